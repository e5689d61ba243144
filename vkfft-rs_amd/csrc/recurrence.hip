// recurrence.hip -- the gated recurrence h[t] = a[t] h[t-1] + m[t] x[t] of every
// channel, and its gradients.
//
// With D the gradient of the state after a token,
//   D[t] = dy[t] + a[t+1] D[t+1],  dx = m D,  da = D (h[t-1] - (m = 1 - a ? x : 0))
// and dgate = da a (1 - a) or da a.
//
// A decay near 1 is kept as what it is short of 1: rounded to 24 bits itself, a
// memory of n tokens would be off by n 2^-25 of its length.
#include <algorithm>

#include "sequence.hpp"
#include "sequence_device.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

// The smaller of a and 1 - a; negative (-0 too) where that is 1 - a.
template <bool SIGMOID>
__device__ __forceinline__ float gate_of(float g) {
    if constexpr (SIGMOID) {
        const float e = expf(-fabsf(g)), small = e / (1.f + e);
        return g > 0.f ? -small : small;
    } else {
        g = g > 0.f ? 0.f : g;  // a NaN stays one
        return g > -0.6931472f ? g == 0.f ? -0.f : expm1f(g) : expf(g);
    }
}
__device__ __forceinline__ bool slow(float s) { return __float_as_int(s) < 0; }
// a v for the gate s.
__device__ __forceinline__ float decayed(float s, float v) { return fmaf(s, v, slow(s) ? v : 0.f); }
__device__ __forceinline__ float short_of(float s) { return slow(s) ? -s : 1.f - s; }  // 1 - a
// da / dgate
template <bool SIGMOID>
__device__ __forceinline__ float slope(float s, float g) {
    if constexpr (SIGMOID) return fabsf(s) * (1.f - fabsf(s));
    return g > 0.f ? 0.f : decayed(s, 1.f);
}

__device__ __forceinline__ long long length(const RecurrenceArgs& a, int b) {
    const long long n = a.lengths ? a.lengths[b] : a.tokens;
    return n < 0 ? 0 : n < a.tokens ? n : a.tokens;
}

template <typename T, bool SIGMOID, bool COMPLEMENT>
__global__ __launch_bounds__(256) void k_recurrence(const RecurrenceArgs a) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    const int b = blockIdx.y;
    if (c >= a.channels) return;
    const long long n = length(a, b), spans = (a.tokens + kSpan - 1) / kSpan;
    const T* x = (const T*)a.x.p + b * a.x.batch + c;
    const T* gate = (const T*)a.gate.p + b * a.gate.batch + c;
    T* y = (T*)a.y.p + b * a.y.batch + c;
    float h = a.state_in ? a.state_in[b * a.channels + c] : 0.f;
    for (long long t = 0; t < a.tokens; ++t) {
        if (a.saved && t % kSpan == 0) a.saved[(b * spans + t / kSpan) * a.channels + c] = h;
        if (t >= n) {
            y[t * a.y.token] = (T)0.f;
            continue;
        }
        const float s = gate_of<SIGMOID>((float)gate[t * a.gate.token]), v = (float)x[t * a.x.token];
        h = decayed(s, h) + (COMPLEMENT ? short_of(s) * v : v);
        y[t * a.y.token] = (T)h;
    }
    if (a.state_out) a.state_out[b * a.channels + c] = h;
}

template <typename T, bool SIGMOID, bool COMPLEMENT>
__global__ __launch_bounds__(256) void k_recurrence_back(const RecurrenceArgs a) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    const int b = blockIdx.y;
    if (c >= a.channels) return;
    const long long n = length(a, b), spans = (a.tokens + kSpan - 1) / kSpan;
    const T* x = (const T*)a.x.p + b * a.x.batch + c;
    const T* gate = (const T*)a.gate.p + b * a.gate.batch + c;
    const T* dy = (const T*)a.dy.p + b * a.dy.batch + c;
    T* dx = (T*)a.y.p + b * a.y.batch + c;
    T* dgate = (T*)a.dgate.p + b * a.dgate.batch + c;
    for (long long t = n; t < a.tokens; ++t) dx[t * a.y.token] = dgate[t * a.dgate.token] = (T)0.f;
    float e = a.state_in ? a.state_in[b * a.channels + c] : 0.f;  // gradient that arrives from the tokens behind
    for (long long span = (n + kSpan - 1) / kSpan - 1; span >= 0; --span) {
        const long long t0 = span * kSpan;
        float s[kSpan], before[kSpan], h = a.saved[(b * spans + span) * a.channels + c];
#pragma unroll
        for (int i = 0; i < kSpan; ++i) {
            const long long t = t0 + i < n ? t0 + i : n - 1;
            s[i] = gate_of<SIGMOID>((float)gate[t * a.gate.token]);
            const float v = (float)x[t * a.x.token];
            before[i] = h;
            h = decayed(s[i], h) + (COMPLEMENT ? short_of(s[i]) * v : v);
        }
#pragma unroll
        for (int i = kSpan - 1; i >= 0; --i) {
            const long long t = t0 + i;
            if (t >= n) continue;
            const float d = (float)dy[t * a.dy.token] + e;
            const float v = (float)x[t * a.x.token], g = (float)gate[t * a.gate.token];
            dx[t * a.y.token] = (T)(COMPLEMENT ? short_of(s[i]) * d : d);
            dgate[t * a.dgate.token] = (T)(d * (COMPLEMENT ? before[i] - v : before[i]) * slope<SIGMOID>(s[i], g));
            e = decayed(s[i], d);
        }
    }
    if (a.state_out) a.state_out[b * a.channels + c] = e;
}

template <typename T, bool SIGMOID, bool COMPLEMENT>
int launch_as(const RecurrenceArgs& a, hipStream_t s, bool back) {
    const auto kernel = back ? k_recurrence_back<T, SIGMOID, COMPLEMENT> : k_recurrence<T, SIGMOID, COMPLEMENT>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.channels + 255) / 256), (unsigned)a.batch), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

template <typename T>
int pick(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.gate_kind == VKFX_GATE_SIGMOID) return a.complement ? launch_as<T, true, true>(a, s, back) : launch_as<T, true, false>(a, s, back);
    return a.complement ? launch_as<T, false, true>(a, s, back) : launch_as<T, false, false>(a, s, back);
}

int pick_element(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return pick<float>(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return pick<_Float16>(a, s, back);
    return pick<__bf16>(a, s, back);
}

}  // namespace

int launch_recurrence_forward(const RecurrenceArgs& a, hipStream_t s) { return pick_element(a, s, false); }
int launch_recurrence_backward(const RecurrenceArgs& a, hipStream_t s) { return pick_element(a, s, true); }
size_t recurrence_workspace_bytes(int, long long, int) { return 16; }

}  // namespace vkfx
