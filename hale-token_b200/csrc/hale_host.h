// hale_host.h -- what the host sides of the library's translation units share:
// the context, error reporting, launch bookkeeping.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <map>
#include <mutex>
#include <set>
#include <string>
#include <utility>
#include <vector>

#include "../../include/hale_cuda.h"

struct hale_comm;

struct hale_ctx {
    int device = 0;
    // objects made on this context; destroying the context detaches them
    // (their own destroy then frees their memory on their device)
    std::set<hale_matrix*> matrices;
    std::set<hale_pool*> pools;
    std::set<hale_decoder*> decoders;
    std::set<hale_comm*> comms;
    int sm_count = 0;
    // expert kernel family (hale_ctx_set_expert_kernel): HALE_EXPERT_AUTO =
    // by batch shape, _TC = tcgen05 kernels, _DP4A = per-CTA kernels (dp4a /
    // warp MMA), _PS = persistent streaming warp-MMA kernels; each where the
    // shapes allow, else the per-CTA kernels
    int expert_kernel = 0;
    std::string msg;
    hale_status status = HALE_OK;
    uint32_t* d_err = nullptr;
    // MoE / route workspace (capacity-based layout; counters first)
    void* ws = nullptr;
    size_t ws_bytes = 0;
    int capM = 0, capE = 0, capK = 0, capH = 0, capI = 0;
    // scratch for unit-level calls
    void* scratch = nullptr;
    size_t scratch_bytes = 0;
    // workspace of the cache and verification calls (hale_serving.cu): made
    // once at its final size, so captured graphs' addresses stay good
    void* serving_ws = nullptr;
    // bumped whenever ws or scratch is reallocated: CUDA graphs captured
    // before hold the old addresses and must not be replayed
    uint64_t ws_gen = 1;
    // hale_moe_forward_host replays: one captured graph per (pool, layer,
    // M, host buffers), valid while ws_gen matches
    struct HostGraph {
        const hale_pool* pool;
        hale_moe_layer layer;
        uint32_t M;
        const void *x, *out, *idx, *w;
        uint64_t gen;
        cudaGraphExec_t exec;
    };
    std::vector<HostGraph> host_graphs;
    cudaStream_t cap_st = nullptr;
    uint32_t* h_err = nullptr;  // page-locked copy of d_err
    uint64_t launches = 0;
    // per-kernel event timing (hale_ctx_profile)
    bool profiling = false;
    struct Mark {
        std::string name;
        cudaEvent_t a, b;
    };
    std::vector<Mark> marks;
    std::vector<cudaEvent_t> spare;
    std::map<std::string, std::pair<uint64_t, double>> totals;
};

// Records the message and status of a failure (on ctx, if any, and for this
// host thread) and returns the status.
hale_status fail(hale_ctx* ctx, hale_status st, const char* fmt, ...);

#define CUDA_TRY(ctx, call)                                                                    \
    do {                                                                                       \
        cudaError_t e_ = (call);                                                               \
        if (e_ != cudaSuccess)                                                                 \
            return fail((ctx), e_ == cudaErrorMemoryAllocation ? HALE_E_OUT_OF_MEMORY : HALE_E_CUDA, \
                        "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__);  \
    } while (0)

inline hale_status check_launch(hale_ctx* ctx, const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(ctx, HALE_E_CUDA, "launch of %s failed: %s", what, cudaGetErrorString(e));
    ctx->launches++;
    return HALE_OK;
}

inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// Opts a kernel into more than 48 KB of dynamic shared memory (once per
// kernel and size; the attribute is per function, not per launch).
// Static shared memory counts toward the same 48 KB default, so the opt-in
// is made for every dynamic size, cached per device and function.
template <class F>
cudaError_t allow_smem(F* func, size_t bytes) {
    if (bytes == 0) return cudaSuccess;
    static std::mutex mu;
    static std::map<std::pair<int, const void*>, size_t> granted;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    size_t& g = granted[{dev, reinterpret_cast<const void*>(func)}];
    if (bytes <= g) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) g = bytes;
    return e;
}

inline cudaEvent_t take_event(hale_ctx* ctx) {
    if (!ctx->spare.empty()) {
        cudaEvent_t e = ctx->spare.back();
        ctx->spare.pop_back();
        return e;
    }
    cudaEvent_t e = nullptr;
    cudaEventCreate(&e);
    return e;
}

// Brackets one launch with events when profiling is on.
struct ProfScope {
    hale_ctx* ctx;
    const char* name;
    cudaStream_t st;
    cudaEvent_t a = nullptr;
    ProfScope(hale_ctx* c, const char* n, cudaStream_t s) : ctx(c), name(n), st(s) {
        if (ctx->profiling) {
            a = take_event(ctx);
            cudaEventRecord(a, st);
        }
    }
    ~ProfScope() {
        if (a) {
            cudaEvent_t b = take_event(ctx);
            cudaEventRecord(b, st);
            ctx->marks.push_back({name, a, b});
        }
    }
};

inline bool stream_capturing(void* stream) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(S(stream), &cs) != cudaSuccess) return false;
    return cs != cudaStreamCaptureStatusNone;
}

inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
// Dynamic shared memory one CTA may ask for on sm_100 (227 KB).
static constexpr size_t kMaxDynSmem = 227 * 1024;
inline bool is_float(hale_dtype d) { return d == HALE_F32 || d == HALE_F16 || d == HALE_BF16; }
inline int float_code(hale_dtype d) { return d == HALE_F32 ? 0 : (d == HALE_F16 ? 1 : 2); }
