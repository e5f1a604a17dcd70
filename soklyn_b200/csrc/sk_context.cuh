// The context behind the C ABI and what every entry point does with it: error texts, launch timing.
#pragma once

#include <cstdarg>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cuda.h>
#include <cuda_runtime.h>
#include <map>
#include <tuple>
#include <vector>

#include "../../include/soklyn_b200.h"

namespace sk { struct TcSplitMaps; }

struct sk_ctx {
    int device = 0;
    uint32_t tile_dim = 16;
    cudaStream_t stream = nullptr;
    bool own_stream = false;
    void *workspace = nullptr;
    size_t workspace_bytes = 0;
    int num_sms = 148;
    size_t smem_optin = 0;
    uint64_t launches = 0;
    char err[512] = {0};
    // tensor-core path
    int cc_major = 0;
    uint32_t gemm_engine = 0;              // 0 auto, 1 FFMA only
    int *tc_err = nullptr;                 // device word a tcgen05 kernel sets when a bounded wait gives up
    int *loss_err = nullptr;               // the word behind it: bits of the losses' indices out of range
    uint64_t loss_launches = 0;
    void *encode_tiled = nullptr;          // cuTensorMapEncodeTiled, resolved through the runtime
    std::map<std::tuple<const void *, uint64_t, uint64_t, uint64_t, uint32_t, uint32_t>, CUtensorMap> tmaps;
    uint64_t tc_launches = 0;
    uint32_t tc_group_n = 8;               // tile columns walked together (SK_TC_GROUP_N at context creation)
    uint32_t handover_min_rows = 0;        // column sums ride in the dX epilogue from this many rows on (SK_HANDOVER_MIN_ROWS at context creation)
    uint32_t reserve_sms = 0;              // SMs the tensor-core GEMMs leave free (for a concurrent exchange kernel)
    uint32_t cluster_blocks[4] = {0, 0, 0, 0};   // blocks the chip holds at once in clusters of 1, 2, 4, 8 (one block per SM; 0: none)
    bool lean = false;                     // SK_OPTION_LEAN_BACKWARD
    // data-parallel backward
    uint32_t *dp_counters = nullptr;       // one completion counter per (layer, block), zero between launches
    // f32 GEMMs on the tensor cores (SK_OPTION_F32_TENSOR_CORES): device copies of the tensor maps of a launch
    bool f32_tensor = false;
    sk::TcSplitMaps *split_maps = nullptr; // ring of kSplitMapSlots entries
    uint32_t split_slot = 0;
    // Column sums handed from the dX epilogue to the weight update of the same layer. Only inside
    // sk_ffn_backward (nothing can touch the tensors or the workspace in between there).
    bool in_ffn_backward = false;
    bool colsum_handover = false;             // SK_OPTION_COLSUM_HANDOVER
    const void *fused_colsum_key = nullptr;   // d_prenorm of the layer whose partial sums sit in the workspace
    uint32_t fused_colsum_groups = 0, fused_colsum_batch = 0;
    // whole-step graphs (sk_step_begin / sk_step_end)
    struct StepGraph { cudaGraphExec_t exec = nullptr; bool warmed = false; uint64_t shape = 0; };   // shape: launch_shape of the record
    StepGraph step_graphs[SK_STEP_SLOTS];
    int step_open = -1;                    // slot between begin and end
    bool step_capturing = false;
    bool allocating = false;               // between sk_step_allocations(1) and (0), with the capture mode the thread had
    cudaStreamCaptureMode caller_mode = cudaStreamCaptureModeGlobal;
    cudaStream_t record_stream = nullptr;  // the calls of a step are recorded on this stream (the legacy default stream
    cudaStream_t user_stream = nullptr;    // cannot be captured); `stream` points here meanwhile, user_stream keeps the caller's
    uint64_t step_stats[4] = {0, 0, 0, 0}; // instantiated, updated in place, launched, unrecorded steps
    // optional per-class event timing
    bool profiling = false;
    std::vector<cudaEvent_t> ev_pool;      // pairs: [2i] start, [2i+1] stop
    std::vector<uint32_t> ev_class;        // class of pair i
    size_t ev_used = 0;
};

namespace sk {

inline int fail(sk_ctx *c, int code, const char *fmt, ...) {
    if (c) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(c->err, sizeof c->err, fmt, ap);
        va_end(ap);
    }
    return code;
}

inline int step_recording(sk_ctx *c) {
    return fail(c, SK_ERR_INVALID_CONFIGURATION, "not while a step graph is being recorded (sk_step_end or sk_step_abort first)");
}

inline int check_cuda(sk_ctx *c, cudaError_t e, const char *what) {
    if (e == cudaSuccess) return SK_OK;
    return fail(c, SK_ERR_DRIVER, "%s: %s", what, cudaGetErrorString(e));
}

// Brackets one launch with events when profiling is on.
struct ProfScope {
    sk_ctx *c;
    size_t slot = (size_t)-1;
    cudaStream_t st;
    ProfScope(sk_ctx *ctx, uint32_t cls, cudaStream_t on = nullptr) : c(ctx), st(on ? on : ctx->stream) {
        if (!c->profiling) return;
        if (c->ev_used * 2 + 2 > c->ev_pool.size()) {
            cudaEvent_t a, b;
            if (cudaEventCreate(&a) != cudaSuccess || cudaEventCreate(&b) != cudaSuccess) return;
            c->ev_pool.push_back(a); c->ev_pool.push_back(b); c->ev_class.push_back(cls);
        }
        slot = c->ev_used++;
        c->ev_class[slot] = cls;
        cudaEventRecord(c->ev_pool[2 * slot], st);
    }
    ~ProfScope() { if (slot != (size_t)-1) cudaEventRecord(c->ev_pool[2 * slot + 1], st); }
};

} // namespace sk
