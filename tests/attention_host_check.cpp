// The host side of the attention operators (vw_api.cpp, vw_attention.cpp) over a CUDA runtime and kernels that only keep
// a record: which memory a launch was given, what was freed, cleared, waited for and recorded, and in which order.
// Compiled and run by tests/test_attention_host.py; argv[1] names a scenario, the exit status says whether it held.

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <set>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "vwsampler.h"
#include "vw_attention.h"
#include "vw_handle.h"
#include "vw_internal.h"

// ------------------------------------------------------------------------------------------------ the recording runtime
struct Op {
    std::string what;        // "malloc", "free", "memset", "device sync", "stream sync", "wait", "record", "launch"
    cudaStream_t stream;
    const void* ptr;         // memory, or the event
    size_t bytes;
};
static std::vector<Op> ops;
static std::map<char*, size_t> live;                 // device memory
static std::map<char*, size_t> freed;
static std::set<void*> pinned;
static std::set<const void*> upload_sources;         // pinned memory that a captured copy reads
static std::set<cudaStream_t> capturing;
static std::set<cudaEvent_t> recorded;
static uintptr_t next_handle = 0x1000;
static unsigned* late_word = nullptr;                // gets late_bits when the host next waits for a stream
static unsigned late_bits = 0;
static cudaError_t next_launch = cudaSuccess;        // what the next decode launch returns

static void note(const char* what, cudaStream_t st = nullptr, const void* p = nullptr, size_t n = 0) {
    ops.push_back({what, st, p, n});
}
static size_t count(const char* what, size_t from = 0) {
    size_t n = 0;
    for (size_t i = from; i < ops.size(); ++i) n += ops[i].what == what;
    return n;
}
static cudaStreamCaptureMode mode = cudaStreamCaptureModeGlobal;
static cudaError_t unless_capturing() {
    return capturing.empty() || mode == cudaStreamCaptureModeRelaxed ? cudaSuccess : cudaErrorStreamCaptureUnsupported;
}

extern "C" {
cudaError_t cudaGetDeviceCount(int* n) { return *n = 1, cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { return *v = 0, cudaSuccess; }
cudaError_t cudaGetDeviceProperties(cudaDeviceProp* p, int) {
    std::memset(p, 0, sizeof *p);
    p->major = 10;
    p->multiProcessorCount = 148;
    return cudaSuccess;
}
const char* cudaGetErrorString(cudaError_t) { return "recorded error"; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes*, const void*) { return cudaErrorInvalidValue; }
cudaError_t cudaMalloc(void** p, size_t n) {
    if (unless_capturing() != cudaSuccess) return cudaErrorStreamCaptureUnsupported;
    *p = std::calloc(n, 1);
    live[static_cast<char*>(*p)] = n;
    note("malloc", nullptr, *p, n);
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
    if (!p) return cudaSuccess;
    auto it = live.find(static_cast<char*>(p));
    if (it == live.end()) return cudaErrorInvalidValue;
    freed.insert(*it);   // (kept, so that its address is not given out again)
    live.erase(it);
    note("free", nullptr, p);
    return cudaSuccess;
}
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) {
    if (unless_capturing() != cudaSuccess) return cudaErrorStreamCaptureUnsupported;
    pinned.insert(*p = std::calloc(n, 1));
    return cudaSuccess;
}
cudaError_t cudaMallocHost(void** p, size_t n) { return cudaHostAlloc(p, n, 0); }
cudaError_t cudaFreeHost(void* p) { return pinned.erase(p) ? cudaSuccess : cudaErrorInvalidValue; }   // (kept too)
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { return std::memcpy(d, s, n), cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t st) {
    if (capturing.count(st)) upload_sources.insert(s);
    return std::memcpy(d, s, n), cudaSuccess;
}
cudaError_t cudaMemcpy2DAsync(void*, size_t, const void*, size_t, size_t, size_t, cudaMemcpyKind, cudaStream_t) {
    return cudaSuccess;
}
cudaError_t cudaMemset(void* p, int v, size_t n) { return std::memset(p, v, n), note("memset", nullptr, p, n), cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t st) {
    return std::memset(p, v, n), note("memset", st, p, n), cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() { return note("device sync"), unless_capturing(); }
cudaError_t cudaStreamSynchronize(cudaStream_t st) {
    if (late_word) *late_word |= late_bits;
    late_word = nullptr;
    return note("stream sync", st), unless_capturing();
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) {
    return *s = reinterpret_cast<cudaStream_t>(next_handle += 16), cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus* c) {
    return *c = capturing.count(s) ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone, cudaSuccess;
}
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { return std::swap(*m, mode), cudaSuccess; }
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) { return note("wait", s, e), cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) {
    return *e = reinterpret_cast<cudaEvent_t>(next_handle += 16), cudaSuccess;
}
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { return recorded.insert(e), note("record", s, e), cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
}

// ------------------------------------------------------------------------------------------------- the recording kernels
namespace vw {
static cudaError_t launched(cudaStream_t st, std::initializer_list<const void*> memory) {
    note("launch", st);
    for (const void* p : memory) note("used", st, p);
    return cudaSuccess;
}
cudaError_t launch_apply_penalty(float*, int, const int32_t*, int64_t, float, unsigned*, cudaStream_t st) {
    return launched(st, {});
}
cudaError_t launch_batch_code_embedding(const BatchDevice&, int, const EmbedOut&, unsigned*, cudaStream_t st) {
    return launched(st, {});
}
cudaError_t launch_batch_commit(const BatchDevice&, const int32_t*, int32_t*, const EmbedOut*, unsigned*, cudaStream_t st) {
    return launched(st, {});
}
cudaError_t launch_batch_draw(const BatchDevice&, int, const DevOptions* opts, int, double*, cudaStream_t st) {
    return launched(st, {opts});
}
cudaError_t launch_batch_record_codes(const BatchDevice&, const int32_t*, int, const EmbedOut*, unsigned*, cudaStream_t st) {
    return launched(st, {});
}
cudaError_t launch_exp_diagnostic(const double*, int64_t, double*, double*, int, cudaStream_t st) { return launched(st, {}); }
cudaError_t launch_frame_embedding(const int32_t*, int, int, int, const uint16_t* const*, int, int, const float*, float*,
                                   unsigned*, cudaStream_t st) {
    return launched(st, {});
}
cudaError_t launch_head_gemm(const void*, int64_t, const void*, int64_t, int, int, int, float* out, int64_t, unsigned*,
                             cudaStream_t st) {
    return launched(st, {out});
}
cudaError_t launch_sampler(const LaunchParams& p, const LaunchPlan&, cudaStream_t st) {
    return launched(st, {p.gscratch, p.deferred_rows, p.deferred_count, p.dev_opts});
}
bool plan_launch(LaunchParams&, int, int, LaunchPlan* plan) {
    *plan = LaunchPlan{8, 8, 1024, 1024};
    return true;
}
int64_t sampler_gscratch_stride(int vmax) { return 28 * vmax; }
cudaError_t static_scratch_address(char**) { return cudaErrorInvalidValue; }
cudaError_t clear_error_bits(unsigned* err, unsigned bits, cudaStream_t st) {
    *err &= ~bits;
    note("clear bits", st, err, bits);
    return cudaSuccess;
}

// sizes that follow the call's, as the kernels' own plans do
TilePlan plan_prompt(const AttnParams& a, int sms) {
    return {1, sms, 128, int64_t{a.batch.n_rows} * a.rows.n_q_heads + 256 * sms, a.batch.n_seqs};
}
TilePlan plan_prefix(const AttnParams& a, int sms) {
    return {1, sms, 128, int64_t{a.batch.n_seqs} * a.rows.n_q_heads + 256 * sms, a.prefix.n_groups};
}
DecodePlan plan_decode(const AttnParams& a, int sms) {
    const int64_t items = int64_t{a.batch.n_seqs} * a.cache.n_kv_heads;
    return {2 * sms, sms, 2, 1, 128, items, (items + 2 * sms) * 2};
}
static cudaError_t tiles(const TileWork& w, cudaStream_t st) {
    return launched(st, {w.counters, w.units_per_cta, w.unit_end, w.part_lse, w.part_o});
}
cudaError_t launch_prompt_attention(const AttnParams&, const TilePlan&, const TileWork& w, cudaStream_t st) {
    return tiles(w, st);
}
cudaError_t launch_prefix_attention(const AttnParams&, const TilePlan&, const TileWork& w, cudaStream_t st) {
    return tiles(w, st);
}
cudaError_t launch_decode_attention(const AttnParams&, const DecodePlan&, const DecodeWork& w, cudaStream_t st) {
    if (next_launch != cudaSuccess) return next_launch;
    return launched(st, {w.tickets, w.units_per_cta, w.unit_end, w.chunk, w.part_lse, w.part_o});
}
cudaError_t launch_rope_append(const RopeParams&, int, cudaStream_t st) { return launched(st, {}); }
}  // namespace vw

// ------------------------------------------------------------------------------------------------------------- scenarios
static int failures = 0;
static void expect(bool ok, const char* what) {
    if (ok) return;
    std::printf("failed: %s\n", what);
    ++failures;
}
static const void* in_freed(size_t from, size_t to) {   // memory that the launches ops[from, to) were given, freed since
    for (size_t i = from; i < to; ++i)
        if (ops[i].what == "used" && ops[i].ptr)
            for (const auto& f : freed)
                if (ops[i].ptr >= f.first && ops[i].ptr < f.first + f.second) return ops[i].ptr;
    return nullptr;
}

struct Calls {
    vw_handle* h = nullptr;
    alignas(64) char memory[256] = {};   // stands for every tensor: nothing reads it
    Calls() { expect(vw_create(0, &h) == VW_OK, "vw_create"); }
    int32_t* ints() { return reinterpret_cast<int32_t*>(memory); }
    vw_kv_cache cache() { return {memory, memory, 16 * 8 * 128, 8 * 128, 128, 1000, 16, 8, 128}; }
    vw_kv_batch batch(int seqs, int rows) { return {ints(), 100, 100, seqs, ints(), ints(), rows}; }
    vw_attn_rows rows() { return {memory, 16 * 128, 128, 16, 0.1f, memory, 16 * 128, 128, nullptr}; }
    vw_status prompt(int rows_, cudaStream_t st) {
        const vw_kv_cache c = cache();
        const vw_kv_batch b = batch(1, rows_);
        const vw_attn_rows r = rows();
        return vw_prompt_attention(h, &c, &b, &r, st);
    }
    vw_status decode(int seqs, cudaStream_t st, int groups = 0) {
        const vw_kv_cache c = cache();
        const vw_kv_batch b = batch(seqs, seqs);
        const vw_attn_rows r = rows();
        const vw_kv_prefix p{ints(), 100, 100, groups, ints(), ints()};
        return vw_decode_attention(h, &c, &b, &p, &r, st);
    }
    vw_status append(int seqs, cudaStream_t st) {
        const vw_kv_cache c = cache();
        const vw_kv_batch b = batch(seqs, seqs);
        vw_rope_rows r{};
        r.q = r.k = r.v = r.q_out = memory;
        r.n_q_heads = 16;
        r.dtype = VW_BF16;
        return vw_rope_append(h, &c, &b, &r, st);
    }
    vw_segment segment(int n, int vocab) {
        vw_segment s{};
        s.logits = memory;
        s.row_stride = s.vocab = vocab;
        s.n_rows = n;
        s.kind = VW_ROWS_SUB;
        s.uniforms = reinterpret_cast<double*>(memory);
        s.out_ids = ints();
        return s;
    }
    vw_status sample(int n, int vocab, int n_options, cudaStream_t st, float penalty = 1.0f) {
        const std::vector<vw_options> o(n_options, vw_options{1, 50, 1.0f, 0.9f, penalty});
        const vw_segment s = segment(n, vocab);
        return vw_sample(h, &s, 1, o.data(), n_options, VW_MEM_DEVICE, st);
    }
    vw_status head(int n, int vocab, cudaStream_t st) {
        const vw_options o{1, 50, 1.0f, 0.9f, 1.0f};
        const vw_segment s = segment(n, vocab);
        return vw_head_sample(h, memory, 64, 64, memory, 64, &s, &o, 1, nullptr, st);
    }
    cudaStream_t stream() {
        cudaStream_t s;
        cudaStreamCreateWithFlags(&s, 0);
        return s;
    }
};

// A graph holds the addresses that its launches were given: no later call may free them before the handle goes.
static void captured_workspace() {
    Calls c;
    cudaStream_t st = c.stream();
    for (int groups : {0, 3}) expect(c.decode(40, st, groups) == VW_OK, "a step before the capture");
    capturing.insert(st);
    const size_t from = ops.size();
    for (int groups : {0, 3}) expect(c.decode(40, st, groups) == VW_OK, "a captured step");
    const size_t to = ops.size();
    capturing.clear();
    for (int rows : {2000, 20000, 100000}) expect(c.prompt(rows, st) == VW_OK, "a prompt that needs more");
    expect(c.decode(5000, st, 3) == VW_OK, "a step that needs more tickets");
    expect(!in_freed(from, to), "memory of a captured step was freed");
    vw_destroy(c.h);
    expect(live.empty(), "the handle leaves nothing allocated");
}
// Without a capture an outgrown buffer goes at once.
static void outgrown_workspace() {
    Calls c;
    cudaStream_t st = c.stream();
    for (int rows = 1000; rows < 200000; rows *= 2) expect(c.prompt(rows, st) == VW_OK, "prompt");
    size_t bytes = 0;
    for (const auto& m : live) bytes += m.second;
    expect(bytes < 2 * size_t{128000} * 16 * 130 * 4, "outgrown buffers are kept");
    vw_destroy(c.h);
    expect(live.empty(), "the handle leaves nothing allocated");
}
// A capture cannot grow the workspace: the call says so and touches nothing; the capture and later calls are not harmed.
static void growth_under_capture() {
    Calls c;
    cudaStream_t st = c.stream();
    for (bool warm : {false, true}) {
        if (warm) expect(c.decode(40, st, 2) == VW_OK && c.prompt(100, st) == VW_OK, "calls before the capture");
        capturing.insert(st);
        const size_t from = ops.size();
        expect(c.decode(4000, st, 2) == VW_ERR_INVALID_ARG, "a captured step that must grow is refused");
        expect(std::string(vw_last_error(c.h)).find("captur") != std::string::npos, "the message says why");
        expect(c.prompt(90000, st) == VW_ERR_INVALID_ARG, "a captured prompt that must grow is refused");
        for (const char* what : {"malloc", "free", "device sync", "stream sync", "memset", "launch"})
            expect(count(what, from) == 0, what);
        if (warm) expect(c.decode(40, st, 2) == VW_OK, "one that fits is captured");
        capturing.clear();
    }
    expect(c.decode(4000, st, 2) == VW_OK, "the same call outside");
    vw_destroy(c.h);
    expect(live.empty(), "the handle leaves nothing allocated");
}

// The same for the sampler's buffers: scratch, deferred rows, the head's logits, a batch's logits, options in a table.
static void captured_sampler() {
    Calls c;
    cudaStream_t st = c.stream();
    const vw_options o{1, 50, 1.0f, 0.9f, 1.0f};
    vw_batch* b = nullptr;
    expect(vw_batch_create(c.h, 4000, 64, 10, 3, 0, 0, 0, &b) == VW_OK, "batch");
    const auto group = [&](int vocab) {
        return vw_batch_sub_head_step(b, 1, c.memory, 64, 64, c.memory, 64, vocab, &o, 1, c.ints(), nullptr, st);
    };
    const auto step = [&] {
        return c.head(16, 64, st) == VW_OK && c.sample(8, 64, 1, st) == VW_OK && group(64) == VW_OK;
    };
    expect(step() && c.sample(8, 64, 40, st) == VW_OK, "before the capture");
    capturing.insert(st);
    const size_t from = ops.size();
    expect(step(), "captured");
    expect(c.sample(8, 64, 40, st, 1.5f) == VW_OK, "captured, with a table of options");
    const size_t to = ops.size();
    capturing.clear();
    expect(group(8192) == VW_OK, "more of a batch's logits");
    expect(c.sample(300000, 4096, 100, st) == VW_OK && c.head(5000, 2048, st) == VW_OK, "calls that need more");
    expect(c.sample(8, 64, 40, st, 1.25f) == VW_OK, "a table as long as the captured one");
    expect(!in_freed(from, to), "memory of a captured call was freed");
    for (const void* p : upload_sources) {
        expect(pinned.count(const_cast<void*>(p)) == 1, "the source of a captured upload was freed");
        expect(static_cast<const vw_options*>(p)->repetition_penalty == 1.5f, "the source of a captured upload was overwritten");
    }
    expect(upload_sources.size() == 1, "one captured upload");
    vw_batch_destroy(b);
    vw_destroy(c.h);
    expect(live.empty() && pinned.empty(), "the handle leaves nothing allocated");
}

static size_t clears(const char* base, size_t bytes, size_t from) {   // of memory [base, base + bytes) since ops[from]
    size_t n = 0;
    for (size_t i = from; i < ops.size(); ++i) {
        const char* p = static_cast<const char*>(ops[i].ptr);
        n += ops[i].what == "memset" && p >= base && p < base + bytes;
    }
    return n;
}
// An error of one stream's call, read there, leaves alone what a call that runs on another stream counts with, and an
// error that arrives meanwhile.  Only a wait that gave up leaves counters to clear, once nothing runs.
static void error_on_another_stream() {
    Calls c;
    cudaStream_t a = c.stream(), b = c.stream();
    expect(c.decode(40, b, 2) == VW_OK && c.prompt(300, b) == VW_OK && c.sample(8, 64, 1, b) == VW_OK, "calls on one stream");
    for (unsigned bit = 1; bit <= vw::kErrKvLens; bit *= 2) {
        const size_t from = ops.size();
        *c.h->d_err |= bit;
        late_word = c.h->d_err;
        late_bits = bit == vw::kErrPosition ? vw::kErrCodeRange : vw::kErrPosition;
        expect(vw_synchronize(c.h, a) != VW_OK, "an error is reported");
        const size_t cleared = clears(c.h->attn_counts.p, c.h->attn_counts.bytes, from) +
                               clears(c.h->defer.p, c.h->defer.bytes, from);
        if (bit == vw::kErrTimeout) {
            size_t waited = ops.size();
            for (size_t i = ops.size(); i-- > from;)
                if (ops[i].what == "device sync") waited = i;
            expect(cleared == 2 && clears(c.h->attn_counts.p, c.h->attn_counts.bytes, waited) == 1 &&
                       clears(c.h->defer.p, c.h->defer.bytes, waited) == 1,
                   "counters are cleared once nothing runs");
        } else {
            expect(cleared == 0, "counters of another stream's calls were cleared");
        }
        expect(vw_synchronize(c.h, b) != VW_OK, "an error that arrived meanwhile is reported too");
        expect(vw_synchronize(c.h, b) == VW_OK && *c.h->d_err == 0, "each once");
    }
    vw_destroy(c.h);
}

// A call that returns after its work reports what calls enqueued before it left, too.
static void error_of_an_enqueued_call() {
    Calls c;
    vw_batch* b = nullptr;
    expect(vw_batch_create(c.h, 4, 64, 10, 3, 0, 0, 0, &b) == VW_OK, "batch");
    const vw_options o{1, 50, 1.0f, 0.9f, 1.0f};
    const int32_t ids[1] = {0};
    float row[4] = {};
    float* out = reinterpret_cast<float*>(c.memory);
    const uint16_t* table[1] = {reinterpret_cast<uint16_t*>(c.memory)};
    const std::vector<std::pair<const char*, std::function<vw_status()>>> calls = {
        {"prompt", [&] { return c.prompt(20, nullptr); }},
        {"decode", [&] { return c.decode(5, nullptr); }},
        {"decode with a prefix", [&] { return c.decode(5, nullptr, 2); }},
        {"append", [&] { return c.append(5, nullptr); }},
        {"sample", [&] { return c.sample(8, 64, 1, nullptr); }},
        {"head and sample", [&] { return c.head(8, 64, nullptr); }},
        {"head", [&] { return vw_head_logits(c.h, c.memory, 64, 64, c.memory, 64, 8, 64, out, nullptr); }},
        {"batch head", [&] {
             return vw_batch_sub_head_step(b, 1, c.memory, 64, 64, c.memory, 64, 64, &o, 1, c.ints(), nullptr, nullptr);
         }},
        {"code embedding", [&] { return vw_batch_code_embedding(b, 1, c.memory, 8, 8, out, 8, nullptr); }},
        {"frame embedding", [&] {
             return vw_frame_embedding(c.h, c.ints(), 2, 2, 8, table[0], 8, table, 8, nullptr, out, nullptr);
         }},
        {"penalty", [&] { return vw_apply_repetition_penalty(c.h, row, 4, ids, 1, 1.5f, VW_MEM_HOST); }},
    };
    for (const auto& call : calls) {
        expect(call.second() == VW_OK, call.first);
        *c.h->d_err |= vw::kErrPageRange;
        if (call.second() != VW_ERR_OUT_OF_RANGE) {
            expect(false, "an earlier call's error was lost by");
            std::printf("    %s\n", call.first);
        }
        expect(call.second() == VW_OK, "and is reported once");
    }
    vw_batch_destroy(b);
    vw_destroy(c.h);
}

// Attention calls share the workspace: each waits for the one before it, whatever its stream's handle says (a new stream
// may have a destroyed one's), also where that one stopped half way.
static void workspace_order() {
    Calls c;
    cudaStream_t a = c.stream(), b = c.stream();
    const auto waits_for_the_last = [&](const char* what, const std::function<vw_status()>& call, cudaStream_t st) {
        size_t launch = 0;   // the last launch so far, and the record behind it
        for (size_t i = 0; i < ops.size(); ++i)
            if (ops[i].what == "launch") launch = i;
        const void* event = nullptr;
        for (size_t i = launch; i < ops.size(); ++i)
            if (ops[i].what == "record" && ops[i].stream == ops[launch].stream) event = ops[i].ptr;
        const size_t from = ops.size();
        expect(call() == VW_OK, what);
        bool waited = false, launched_before = false;
        for (size_t i = from; i < ops.size(); ++i) {
            launched_before = launched_before || ops[i].what == "launch";
            waited = waited || (!launched_before && ops[i].what == "wait" && ops[i].stream == st && ops[i].ptr == event);
        }
        expect(event && waited, what);
    };
    expect(c.decode(40, a, 2) == VW_OK && c.prompt(300, a) == VW_OK, "first calls");
    waits_for_the_last("on another stream", [&] { return c.decode(40, b, 2); }, b);
    waits_for_the_last("on a stream with the same handle", [&] { return c.decode(40, b, 2); }, b);
    waits_for_the_last("a prompt on it", [&] { return c.prompt(300, b); }, b);
    waits_for_the_last("on the handle's stream", [&] { return c.prompt(300, nullptr); }, c.h->stream);
    next_launch = cudaErrorInvalidValue;
    expect(c.decode(40, a, 2) == VW_ERR_CUDA, "a call whose second kernel does not start");
    next_launch = cudaSuccess;
    waits_for_the_last("after a call that stopped half way", [&] { return c.decode(40, b); }, b);
    // within a capture no event of uncaptured work is waited for, and none is recorded
    capturing.insert(a);
    const size_t from = ops.size();
    expect(c.decode(40, a, 2) == VW_OK && c.prompt(300, a) == VW_OK, "captured");
    expect(count("wait", from) == 0 && count("record", from) == 0, "captured calls are ordered by their graph");
    capturing.clear();
    vw_destroy(c.h);
}

int main(int argc, char** argv) {
    const std::map<std::string, std::function<void()>> scenarios = {
        {"captured_workspace", captured_workspace},
        {"outgrown_workspace", outgrown_workspace},
        {"growth_under_capture", growth_under_capture},
        {"captured_sampler", captured_sampler},
        {"error_on_another_stream", error_on_another_stream},
        {"error_of_an_enqueued_call", error_of_an_enqueued_call},
        {"workspace_order", workspace_order},
    };
    const auto it = argc > 1 ? scenarios.find(argv[1]) : scenarios.end();
    if (it == scenarios.end()) return 2;
    it->second();
    return failures ? 1 : 0;
}
