// vw_tc.cuh -- what the tcgen05 kernels share (vw_head.cu, vw_prompt.cu): bounded mbarrier waits, shared-memory matrix
// descriptors, TMA loads and tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "vw_attention.h"
#include "vw_internal.h"

namespace vw {

__device__ __forceinline__ uint32_t s32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// true once the phase of `parity` completed; false on timeout (sets `err` and `abort`) or when another role aborted
static __device__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int32_t* abort, unsigned* err) {
    if (try_wait(bar, parity)) return true;
    const uint64_t t0 = now_ns();
    while (!try_wait(bar, parity)) {
        if (*abort) return false;
        if (now_ns() - t0 > kWaitLimitNs) {
            atomicOr(err, kErrTimeout);
            *abort = 1;
            return false;
        }
    }
    return true;
}
// the same for a whole warp: one answer for its 32 lanes
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int32_t* abort, unsigned* err) {
    if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait_bounded(bar, parity, abort, err));
}
// the same without a call (where registers are full, a call would spill them)
__device__ __forceinline__ bool spin_warp(uint32_t bar, uint32_t parity, volatile int32_t* abort, unsigned* err) {
    if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
    const uint64_t t0 = now_ns();
    for (;;) {
        if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
        const bool late = now_ns() - t0 > kWaitLimitNs;
        if (__any_sync(0xffffffffu, late || *abort)) {
            if (late) atomicOr(err, kErrTimeout);
            *abort = 1;
            return false;
        }
    }
}
// teardown flavour: bounded, no error reporting (an abort is already recorded)
static __device__ void drain_wait(uint32_t bar, uint32_t parity) {
    const uint64_t t0 = now_ns();
    while (!try_wait(bar, parity))
        if (now_ns() - t0 > kWaitLimitNs) return;
}

// shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row atoms 1024 bytes apart (SBO), version 1
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {   // relative error 2^-22; -inf gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// (by the lanes with `pred`, so that a warp's other code stays uniform)
__device__ __forceinline__ void arrive_if(bool pred, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
        "r"(pred ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ void mma_commit_if(bool pred, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(pred ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda)
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_fn() {
    static std::once_flag once;
    static EncodeTiledFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// row-major [rows, cols] (row pitch `ld` elements of `esize` bytes) in boxes of box_rows x box_cols (128 bytes wide),
// 128-byte swizzle
inline bool make_map(CUtensorMap* m, CUtensorMapDataType type, size_t esize, const void* base, int rows, int cols, int64_t ld,
              int box_rows, int box_cols) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * esize};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    return fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A cache's keys or values in boxes of 64 dims x min(page_size, max_rows) tokens of one head of one page; dims past
// head_dim read zeros
inline bool make_cache_map(CUtensorMap* m, const KvCacheDev& c, const void* base, int max_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size),
                                static_cast<cuuint64_t>(c.n_kv_heads), static_cast<cuuint64_t>(c.n_pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c.token_stride) * 2, static_cast<cuuint64_t>(c.head_stride) * 2,
                                   static_cast<cuuint64_t>(c.page_stride) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(c.page_size < max_rows ? c.page_size : max_rows), 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, ones,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The query rows in boxes of 64 dims x box_heads heads (0: a whole group's) x box_rows rows
inline bool make_row_map(CUtensorMap* m, const AttnParams& a, int box_rows, int box_heads = 0) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.cache.head_dim), static_cast<cuuint64_t>(a.rows.n_q_heads),
                                static_cast<cuuint64_t>(a.batch.n_rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.rows.q_head) * 2, static_cast<cuuint64_t>(a.rows.q_row) * 2};
    const cuuint32_t heads = box_heads ? box_heads : a.rows.n_q_heads / a.cache.n_kv_heads;
    const cuuint32_t box[3] = {64, heads, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t ones[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(a.rows.q), dims, strides, box, ones,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace vw
