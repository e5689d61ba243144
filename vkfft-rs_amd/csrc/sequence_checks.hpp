// sequence_checks.hpp -- what the entry points of the sequence operators share:
// argument checks, plans' memory and lifetime.
#pragma once

#include <algorithm>
#include <exception>
#include <new>
#include <string>

#include "context.hpp"
#include "overlap.hpp"
#include "vkfx.h"

namespace vkfx {

// Runs an entry point's body: no C++ exception leaves the C ABI.
template <typename F>
inline int guarded(F body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(VKFX_ERR_RESOURCE_LIMIT, "out of host memory");
    } catch (const std::exception& ex) {
        return fail(VKFX_ERR_NATIVE_RUNTIME, ex.what());
    }
}

inline int bad(const std::string& what) { return fail(VKFX_ERR_INVALID_ARGUMENT, what); }

inline bool known_element(int32_t e) { return e >= VKFX_ELEMENT_F32 && e <= VKFX_ELEMENT_BF16; }

inline hipStream_t stream_of(const vkfx_context* ctx, void* stream) {
    if (!stream) return ctx->stream;
    return stream == (void*)hipStreamLegacy ? nullptr : (hipStream_t)stream;
}

inline int allocate(DevBuf& b, size_t bytes) {
    if (!bytes) return VKFX_OK;
    const hipError_t e = hipMalloc(&b.p, bytes);
    if (e != hipSuccess) {
        b.p = nullptr;
        return hip_fail(e, "hipMalloc");
    }
    b.bytes = bytes;
    return VKFX_OK;
}

inline void retain(vkfx_context* ctx) {
    std::lock_guard<std::mutex> lock(ctx->mu);
    ++ctx->plans;
}

// Waits for the device: the plan's calls may still run on any stream.
template <typename P>
inline int destroy(P* plan) {
    if (!plan) return VKFX_OK;
    (void)hipSetDevice(plan->ctx->device);
    (void)hipDeviceSynchronize();
    {
        std::lock_guard<std::mutex> lock(plan->ctx->mu);
        --plan->ctx->plans;
    }
    delete plan;
    return VKFX_OK;
}

// The context's device is the current one within a scope; afterwards the one that was.
struct OnDevice {
    int before = -1, device;
    explicit OnDevice(const vkfx_context* ctx) : device(ctx->device) {
        (void)hipGetDevice(&before);
        if (before != device) (void)hipSetDevice(device);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    ~OnDevice() {
        if (before >= 0 && before != device) (void)hipSetDevice(before);
    }
};

// a * b in *out; false past 2^60, from where on a count of bytes could overflow.
inline bool mul(uint64_t a, uint64_t b, uint64_t* out) { return !__builtin_mul_overflow(a, b, out) && *out < (1ull << 60); }

inline uint64_t bytes_of(int32_t element) { return element == VKFX_ELEMENT_F32 ? 4 : 2; }

inline int check_work(const void* d_work) {
    return (uintptr_t)d_work % 16 ? bad("work must be aligned to 16 bytes") : VKFX_OK;
}

// A tensor of a call, for the check that outputs share no memory with inputs
// nor with each other. No data: nothing.
struct Tensor {
    const char* name;
    Region region;
    bool written;
};

inline Tensor flat(const char* name, const void* p, uint64_t bytes, bool written) {
    Tensor t{name, {}, written};
    t.region.at = (uintptr_t)p;
    t.region.run = p ? bytes : 0;
    return t;
}

inline Tensor rows_of(const char* name, const void* p, uint64_t rows, int64_t stride, uint64_t width, int32_t element, bool written) {
    Tensor t = flat(name, p, width * bytes_of(element), written);
    t.region.axis(0, (uint64_t)stride * bytes_of(element), rows);
    return t;
}

inline Tensor sequence_of(const char* name, const vkfx_sequence& s, uint64_t batch, uint64_t tokens, uint64_t heads, uint64_t dim,
                   int32_t element, bool written) {
    const uint64_t size = bytes_of(element);
    Tensor t = flat(name, s.data, dim * size, written);
    t.region.axis(0, (uint64_t)s.batch_stride * size, batch).axis(1, (uint64_t)s.token_stride * size, tokens);
    t.region.axis(2, (uint64_t)s.head_stride * size, heads);
    return t;
}

// `out` and `in`, `out2` and `in2`: the names of outputs that stand in their input's place.
template <size_t N>
inline int check_apart(const Tensor (&tensors)[N], const char* out = nullptr, const char* in = nullptr,
                       const char* out2 = nullptr, const char* in2 = nullptr) {
    uintptr_t end[N];
    for (size_t i = 0; i < N; ++i) end[i] = tensors[i].region.run ? tensors[i].region.at + tensors[i].region.span() : 0;
    for (size_t i = 0; i < N && tensors[i].written; ++i)  // outputs come first
        for (size_t j = i + 1; j < N; ++j) {
            const Tensor &w = tensors[i], &t = tensors[j];
            if (w.region.at >= end[j] || t.region.at >= end[i] || (w.name == out && t.name == in) ||
                (w.name == out2 && t.name == in2))
                continue;
            if (overlap(w.region, t.region)) return bad(std::string(w.name) + " overlaps " + t.name);
        }
    return VKFX_OK;
}

// Strides of one [batch][token][head][dim] tensor: none negative, every offset
// within 62 bits, and for an output no two elements at one place.
inline int check_sequence(const char* name, const vkfx_sequence& s, uint64_t batch, uint64_t tokens, uint64_t heads, uint64_t dim,
                   bool written) {
    if (!s.data) return bad(std::string("null ") + name);
    struct Axis {
        uint64_t stride, extent;
    } axes[3] = {{(uint64_t)s.batch_stride, batch}, {(uint64_t)s.token_stride, tokens}, {(uint64_t)s.head_stride, heads}};
    if (s.batch_stride < 0 || s.token_stride < 0 || s.head_stride < 0) return bad(std::string(name) + ": negative stride");
    std::sort(axes, axes + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    uint64_t span = dim;
    for (const Axis& x : axes) {
        if (x.extent <= 1) continue;
        if (written && x.stride < span) return bad(std::string(name) + ": an output's elements overlap");
        uint64_t reach;
        if (!mul(x.stride, x.extent - 1, &reach) || (span += reach) >= (1ull << 60))
            return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, std::string(name) + ": strides reach past 2^60 elements");
    }
    return VKFX_OK;
}

}  // namespace vkfx
