// What the attention families share: the run workspace and its fences, the
// geometry checks, caller-memory checks (attention.hip: the fp16 cache;
// attention_q8.hip: the 8-bit cache).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cmath>
#include <mutex>

#include "../../include/rk_npu_attention_f16.h"
#include "runtime.hpp"

namespace hm {

constexpr uint32_t MAGIC_ATTN_WORK = 0x57414841u;

// Partial rows a workspace holds: when it splits the keys, plan_attention
// launches fewer than 512 blocks of 64 or 128 query rows, or 1024 of 32 or 4
// (head_dim 256: 64 rows at most).
inline size_t attn_partial_rows(int head_dim) { return (size_t)2048 * (head_dim <= 128 ? 64 : 16); }

// Device-path work (rk_npu_hip_attention_cache_append / _run, enqueued on the
// caller's streams) that a later host call on the same cache or workspace must
// wait for. The host call waits for events after that work, not for the whole
// device:
// - work on the null stream: the event is recorded by the first wait after it.
//   An event costs 4.3 us of the stream's time (its cache flush and signal), a
//   decode step noted three, 25.8 -> 13.6 us without them, and the null stream
//   exists until the process ends and is never captured, so it can be recorded
//   on at any later time;
// - work on another stream, which its owner may destroy or capture afterwards:
//   recorded at once. Work from a second such stream while the first's is still
//   pending, or work under graph capture (whose replays the host cannot see),
//   makes the next wait a device-wide synchronize instead.
struct DevFence {
    std::mutex mu;
    hipEvent_t ev = nullptr;
    hipEvent_t null_ev = nullptr;
    hipStream_t last = nullptr;
    bool used = false;       // ev holds the last work of a stream other than the null stream
    bool null_used = false;  // null_ev holds the null stream's work up to the last wait
    bool null_new = false;   // there is null-stream work since
    bool broad = false;      // wait for the whole device next time

    static bool create(hipEvent_t& e) {
        if (!e && hipEventCreateWithFlags(&e, hipEventDisableTiming) != hipSuccess) {
            (void)hipGetLastError();
            e = nullptr;
        }
        return e != nullptr;
    }
    static bool record(hipEvent_t e, hipStream_t s) {
        if (hipEventRecord(e, s) == hipSuccess) return true;
        (void)hipGetLastError();
        return false;
    }
    // Note device-path work just enqueued on stream s.
    void note(hipStream_t s) {
        std::lock_guard<std::mutex> lock(mu);
        if (!s) {
            null_new = true;
            return;
        }
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone) {
            (void)hipGetLastError();
            broad = true;
            return;
        }
        if (used && s != last) {
            const hipError_t q = hipEventQuery(ev);
            (void)hipGetLastError();  // (not-ready is an answer, not an error)
            if (q != hipSuccess) broad = true;
        }
        if (!create(ev) || !record(ev, s)) {
            broad = true;
            return;
        }
        used = true;
        last = s;
    }
    // Order stream s after the noted work (s == nullptr: the host waits).
    hipError_t wait(hipStream_t s) {
        std::lock_guard<std::mutex> lock(mu);
        if (null_new && !broad) {
            if (create(null_ev) && record(null_ev, nullptr)) {
                null_used = true;
                null_new = false;
            } else {
                broad = true;
            }
        }
        if (broad) {
            const hipError_t e = hipDeviceSynchronize();
            if (e == hipSuccess) broad = used = null_used = null_new = false;
            return e;
        }
        hipError_t e = hipSuccess;
        if (used) e = s ? hipStreamWaitEvent(s, ev, 0) : hipEventSynchronize(ev);
        if (e == hipSuccess && null_used) e = s ? hipStreamWaitEvent(s, null_ev, 0) : hipEventSynchronize(null_ev);
        return e;
    }
    void destroy() {
        if (ev) (void)hipEventDestroy(ev);
        if (null_ev) (void)hipEventDestroy(null_ev);
        ev = null_ev = nullptr;
    }
};

struct AttnWork {
    uint32_t magic;
    Domain* domain;
    rk_npu_attention_f16_config cfg;
    __half* q;     // host-call staging [qh][max_query_rows][D]
    float* out;    // host-call staging (f32; fp16 output uses the first half)
    float* part;   // split partials
    size_t q_bytes, out_bytes, part_bytes;
    hipStream_t stream;
    std::atomic<bool> busy;
    DevFence fence;  // device-path runs writing this workspace's partials
    HostStage hs;    // pinned staging of host-buffer runs
};

// The reference's checks (src/npu.rs:714-728) plus this library's limits.
inline bool valid_config(const rk_npu_attention_f16_config* c) {
    if (!c) return false;
    const int d = c->head_dim;
    return c->kv_heads >= 1 && c->kv_heads <= 32 && c->query_heads >= c->kv_heads &&
           c->query_heads % c->kv_heads == 0 && c->query_heads <= 256 && d > 0 && d % 32 == 0 && d <= 256 &&
           std::isfinite(c->softmax_scale) && c->softmax_scale > 0.0f && c->max_query_rows >= 1 &&
           c->max_query_rows <= 256 && c->max_capacity >= 1 && c->initial_capacity >= 0 &&
           c->initial_capacity <= c->max_capacity &&
           (c->mask_mode == RK_NPU_ATTENTION_F16_CAUSAL || c->mask_mode == RK_NPU_ATTENTION_F16_NO_MASK);
}

// Head dims with a kernel instantiation.
inline bool supported_dim(int d) { return d == 64 || d == 128 || d == 256; }

inline AttnWork* as_attn_work(void* p) {
    AttnWork* w = static_cast<AttnWork*>(p);
    return (w && w->magic == MAGIC_ATTN_WORK) ? w : nullptr;
}

// Whether a kernel on `device` may read caller memory at p: that GPU's own.
// Another GPU's (readable only where peer access is on), managed and host
// memory (pageable memory faults a kernel) keep the copies, which the runtime
// checks and stages.
inline bool kernel_readable(const void* p, int device) {
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return a.type == hipMemoryTypeDevice && a.device == device;
}

}  // namespace hm
