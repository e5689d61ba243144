// context.hpp -- what the C ABI's translation units share: the context, the
// thread's last error and an owned device allocation.
#pragma once

#include <hip/hip_runtime.h>

#include <mutex>
#include <string>
#include <vector>

#include "vkfx.h"

namespace vkfx {

// Message of the last failing call on this thread (vkfx_last_error).
std::string& last_error();

inline int fail(int code, const std::string& msg) {
    last_error() = msg;
    return code;
}

inline int hip_fail(hipError_t e, const char* what) {
    return fail(VKFX_ERR_NATIVE_RUNTIME, std::string(what) + ": " + hipGetErrorString(e));
}

struct DevBuf {
    void* p = nullptr;
    size_t bytes = 0;
    DevBuf() = default;
    DevBuf(const DevBuf&) = delete;
    DevBuf& operator=(const DevBuf&) = delete;
    ~DevBuf() {
        if (p) (void)hipFree(p);
    }
};

}  // namespace vkfx

// Pooled device / pinned host buffer. `ready` (optional) is recorded on the
// stream of its last user; the next user's stream waits on it, so reuse is
// stream-ordered.
struct PoolBuf {
    void* p = nullptr;
    size_t bytes = 0;
    hipEvent_t ready = nullptr;
};

struct vkfx_context {
    int device = 0;
    hipStream_t stream = nullptr;
    vkfx_device_profile profile{};
    std::vector<PoolBuf> dev_pool, host_pool;  // free buffers
    std::vector<hipStream_t> stream_pool;      // free streams for tickets
    void* scratch = nullptr;                   // this device's static scratch (vkfx_execute_noalloc)
    hipError_t scratch_err = hipSuccess;       // why `scratch` is null, if it is
    std::mutex mu;                             // guards the pools, `active` and `plans`
    int active = 0;                            // tickets submitted and not yet destroyed
    int plans = 0;                             // plans (of every kind) created and not yet destroyed
};
