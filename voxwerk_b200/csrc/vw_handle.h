// vw_handle.h -- the handle behind the C ABI and the helpers its entry points share (vw_api.cpp, vw_attention.cpp).
// Not part of the public ABI.
#pragma once

#include <cstddef>
#include <cstdint>
#include <new>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "../../include/vwsampler.h"
#include "vw_internal.h"

#define VW_EXPORT extern "C" __attribute__((visibility("default")))

constexpr int kCopyStreams = 3;   // host -> device copies of VW_MEM_HOST calls run on this many copy engines

// Device memory that grows with a handle's calls.  The kernels of a captured call keep its address for as long as their
// graph lives, so a buffer that a capture has used is put aside when it is outgrown, and freed with the handle.
struct DeviceBuffer {
    char* p = nullptr;
    size_t bytes = 0;
    bool captured = false;
};

struct vw_handle {
    int device = -1;
    cudaStream_t stream = nullptr;
    cudaStream_t copy_streams[kCopyStreams] = {};
    cudaEvent_t copy_events[kCopyStreams + 1] = {};   // one per copy stream, and the fork point
    int sm_count = 0;
    unsigned* d_err = nullptr;      // device error word (kErr* bits)
    unsigned* h_err = nullptr;      // pinned mirror
    DeviceBuffer scratch;           // general-path scratch, one slice per CTA
    DeviceBuffer stage;             // VW_MEM_HOST: device copies of the caller's arrays
    DeviceBuffer logits;            // vw_head_sample: the GEMM's logits when the caller keeps none
    DeviceBuffer defer;             // four counters + the rows the warp-per-row kernel defers
    std::vector<DeviceBuffer> old_defers;   // outgrown ones that captured calls still use
    vw::DevOptions* d_opts = nullptr;
    vw::DevOptions* h_opts = nullptr;   // pinned upload buffer for option tables > kInlineOptions
    std::vector<vw::DevOptions*> captured_opts;   // upload buffers of captured calls, one each
    size_t opts_cap = 0;
    cudaEvent_t opts_done = nullptr;
    unsigned long long* d_stats = nullptr;   // vw::kNumStats per-path row counters
    unsigned long long* d_guess = nullptr;   // candidate thresholds carried from call to call
    int force_exact = 0;                     // VW_FORCE_EXACT at creation
    int test_stall_row = -1;                 // VW_TEST_STALL_ROW at creation (first vw_sample call only)
    unsigned long long h2d_bytes = 0;        // host -> device input bytes of VW_MEM_HOST calls (vw_stats.h2d_bytes)
    DeviceBuffer attn;                       // attention: partial results (vw_attention.cpp)
    DeviceBuffer attn_counts;                // attention: counters and tickets, zero between calls
    std::vector<DeviceBuffer> old_attn_counts;   // outgrown ones that captured calls still use
    std::vector<DeviceBuffer> old_buffers;       // likewise, of any other use
    cudaEvent_t attn_done = nullptr;         // the end of the last call that used them
    std::vector<vw_batch*> batches;          // live batches created on this handle (released by vw_destroy)
    std::string last_error;
};

// Restores the caller's current device on scope exit.
class DeviceGuard {
  public:
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
        if (prev_ == dev) {   // nothing to set or to restore
            prev_ = -1;
            ok_ = true;
            return;
        }
        ok_ = cudaSetDevice(dev) == cudaSuccess;
    }
    ~DeviceGuard() {
        if (prev_ >= 0) cudaSetDevice(prev_);
    }
    bool ok() const { return ok_; }

  private:
    int prev_ = -1;
    bool ok_ = false;
};

inline vw_status fail(vw_handle* h, vw_status s, const std::string& msg) {
    if (h) h->last_error = msg;
    return s;
}

inline vw_status cuda_fail(vw_handle* h, cudaError_t e, const char* where) {
    return fail(h, VW_ERR_CUDA, std::string(where) + ": " + cudaGetErrorString(e));
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

inline size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Lets an outgrown buffer go: put aside where captured calls use it, else freed (the caller has waited for its users).
inline vw_status let_go(vw_handle* h, DeviceBuffer* b, std::vector<DeviceBuffer>* aside, const char* what) {
    if (!b->p) return VW_OK;
    if (b->captured) {
        try {
            aside->push_back(*b);
        } catch (const std::bad_alloc&) {
            return fail(h, VW_ERR_CUDA, what);
        }
    } else {
        const cudaError_t e = cudaFree(b->p);
        if (e != cudaSuccess) return cuda_fail(h, e, what);
    }
    *b = DeviceBuffer{};
    return VW_OK;
}

// Whether work enqueued on `st` goes into a CUDA graph instead of running.
inline bool is_capturing(cudaStream_t st) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(st, &cap) == cudaSuccess && cap != cudaStreamCaptureStatusNone;
}

// Grows a buffer of the handle to `need` bytes, for a call that is being captured or not.  The old one is freed when the
// device is done with it; inside a capture, where that cannot be waited for, it is put aside.
inline vw_status grow(vw_handle* h, DeviceBuffer* b, size_t need, const char* what, bool capturing = false,
                      std::vector<DeviceBuffer>* aside = nullptr) {
    if (need <= b->bytes) {
        b->captured = b->captured || capturing;
        return VW_OK;
    }
    if (b->p) {
        b->captured = b->captured || capturing;
        const cudaError_t e = capturing ? cudaSuccess : cudaDeviceSynchronize();
        if (e != cudaSuccess) return cuda_fail(h, e, what);
        const vw_status r = let_go(h, b, aside ? aside : &h->old_buffers, what);
        if (r != VW_OK) return r;
    }
    const size_t n = round_up(need + need / 4, 1 << 20);
    const cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&b->p), n);
    if (e != cudaSuccess) return cuda_fail(h, e, what);
    b->bytes = n;
    b->captured = capturing;
    return VW_OK;
}

// Waits for `st` and turns, then clears, the device error word.
vw_status read_device_error(vw_handle* h, cudaStream_t st);
