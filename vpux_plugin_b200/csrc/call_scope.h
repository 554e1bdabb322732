// What every entry point that enqueues work does around it: the context's lock and device, the error flags, the
// launch statistics, and the choice between waiting and returning with the work still in flight.
#pragma once

#include <cstring>
#include <mutex>

#include "common.h"

namespace vf {

struct CallScope {  // per-call bookkeeping: context lock, device, error flags, launch statistics
    vf_ctx* ctx;
    std::unique_lock<std::mutex> lock;
    DeviceGuard dev;
    uint64_t launches0;
    vf_stats* stats;
    CallScope(vf_ctx* c, vf_stats* s): ctx(check(c)), lock(c->mu), dev(c->device), launches0(c->launches), stats(s) {
        if (stats) std::memset(stats, 0, sizeof(*stats));
        flags_begin(ctx);
        if (stats && ctx->time_ev[0]) cudaEventRecord(ctx->time_ev[0], ctx->stream);
    }
    static vf_ctx* check(vf_ctx* c) {
        if (!c) raise(VF_ERR_INVALID_ARG, "ctx is NULL");
        return c;
    }
    bool finished = false;
    bool may_defer = false;  // set by calls that touched device memory only
    void finish() {
        if (may_defer && (ctx->opt_flags & VF_OPT_ASYNC)) {
            VF_CUDA(cudaGetLastError());
            ctx->deferred = true;  // the next synchronising call reports what these kernels found
        } else {
            const bool timed = stats && ctx->time_ev[0] && ctx->stream == ctx->main_stream;
            if (timed) cudaEventRecord(ctx->time_ev[1], ctx->stream);
            flags_check(ctx);
            if (timed) cudaEventElapsedTime(&stats->device_ms, ctx->time_ev[0], ctx->time_ev[1]);
        }
        finished = true;
        if (stats) stats->kernels_launched = int32_t(ctx->launches - launches0);
    }
    // A call that ends early (an exception on its way to the caller) still waits for what it enqueued: the
    // caller's buffers and the context's job-table area must not be in use once the call has returned. While the stream is
    // recorded into a graph nothing of it runs, and a wait would end the recording.
    ~CallScope() {
        if (finished) return;
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(ctx->main_stream, &capture) != cudaSuccess || capture != cudaStreamCaptureStatusNone) {
            cudaGetLastError();
            return;
        }
        cudaStreamSynchronize(ctx->main_stream);
        if (ctx->lane_stream) cudaStreamSynchronize(ctx->lane_stream);
        if (ctx->launches != launches0) flags_drop(ctx);
        cudaGetLastError();
    }
};

}  // namespace vf
