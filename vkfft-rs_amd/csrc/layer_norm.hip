// layer_norm.hip -- layer norm of rows and its gradients.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "sequence.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float block_sum(float v, float* lds) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void k_norm_forward(const NormArgs a) {
    __shared__ float lds[4];
    const long long r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.x_stride;
    T* y = (T*)a.y + r * a.y_stride;
    float s = 0.f;
    for (int i = threadIdx.x; i < a.width; i += 256) s += to_f32(x[i]);
    const float mean = block_sum(s, lds) / (float)a.width;
    s = 0.f;
    for (int i = threadIdx.x; i < a.width; i += 256) {
        const float d = to_f32(x[i]) - mean;
        s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, lds) / (float)a.width + a.epsilon);
    for (int i = threadIdx.x; i < a.width; i += 256) {
        const float w = a.weight ? to_f32(((const W*)a.weight)[i]) : 1.f;
        const float b = a.bias ? to_f32(((const W*)a.bias)[i]) : 0.f;
        y[i] = (T)((to_f32(x[i]) - mean) * rstd * w + b);
    }
    if (a.stats_out && threadIdx.x == 0) {
        a.stats_out[2 * r] = mean;
        a.stats_out[2 * r + 1] = rstd;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void k_norm_backward_x(const NormArgs a) {
    __shared__ float lds[4];
    const long long r = blockIdx.x;
    const T* x = (const T*)a.x + r * a.x_stride;
    const T* dy = (const T*)a.dy + r * a.dy_stride;
    T* dx = (T*)a.y + r * a.y_stride;
    const float mean = a.stats_in[2 * r], rstd = a.stats_in[2 * r + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < a.width; i += 256) {
        const float g = to_f32(dy[i]) * (a.weight ? to_f32(((const W*)a.weight)[i]) : 1.f);
        s1 += g;
        s2 += g * ((to_f32(x[i]) - mean) * rstd);
    }
    s1 = block_sum(s1, lds) / (float)a.width;
    s2 = block_sum(s2, lds) / (float)a.width;
    for (int i = threadIdx.x; i < a.width; i += 256) {
        const float g = to_f32(dy[i]) * (a.weight ? to_f32(((const W*)a.weight)[i]) : 1.f);
        dx[i] = (T)((g - s1 - (to_f32(x[i]) - mean) * rstd * s2) * rstd);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_backward_rows(const NormArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    float dw = 0.f, db = 0.f;
    for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float g = to_f32(((const T*)a.dy)[r * a.dy_stride + c]);
        dw += g * (to_f32(((const T*)a.x)[r * a.x_stride + c]) - a.stats_in[2 * r]) * a.stats_in[2 * r + 1];
        db += g;
    }
    a.partial[(long long)blockIdx.y * 2 * a.width + c] = dw;
    a.partial[((long long)blockIdx.y * 2 + 1) * a.width + c] = db;
}

template <typename W>
__global__ __launch_bounds__(256) void k_norm_backward_sum(const NormArgs a, int parts) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    float dw = 0.f, db = 0.f;
    for (int p = 0; p < parts; ++p) {
        dw += a.partial[(long long)p * 2 * a.width + c];
        db += a.partial[((long long)p * 2 + 1) * a.width + c];
    }
    if (a.dweight) ((W*)a.dweight)[c] = (W)dw;
    if (a.dbias) ((W*)a.dbias)[c] = (W)db;
}

constexpr int kParts = 64;

template <typename T, typename W>
int forward_as(const NormArgs& a, hipStream_t s) {
    if (a.rows) hipLaunchKernelGGL((k_norm_forward<T, W>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

template <typename T, typename W>
int backward_as(const NormArgs& a, hipStream_t s) {
    // dx may overwrite dy: the sums over the rows go first
    if (a.dweight || a.dbias) {
        const unsigned cols = (unsigned)((a.width + 255) / 256);
        const int parts = (int)(a.rows < kParts ? a.rows : kParts);
        if (parts) hipLaunchKernelGGL((k_norm_backward_rows<T>), dim3(cols, parts), dim3(256), 0, s, a);
        hipLaunchKernelGGL((k_norm_backward_sum<W>), dim3(cols), dim3(256), 0, s, a, parts);
    }
    if (a.y && a.rows) hipLaunchKernelGGL((k_norm_backward_x<T, W>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

template <typename T>
int pick(const NormArgs& a, hipStream_t s, bool forward) {
    if (a.weight_element == VKFX_ELEMENT_F32) return forward ? forward_as<T, float>(a, s) : backward_as<T, float>(a, s);
    return forward ? forward_as<T, T>(a, s) : backward_as<T, T>(a, s);
}

int pick_element(const NormArgs& a, hipStream_t s, bool forward) {
    if (a.element == VKFX_ELEMENT_F32) return pick<float>(a, s, forward);
    if (a.element == VKFX_ELEMENT_F16) return pick<_Float16>(a, s, forward);
    return pick<__bf16>(a, s, forward);
}

}  // namespace

int launch_norm_forward(const NormArgs& a, hipStream_t s) { return pick_element(a, s, true); }
int launch_norm_backward(const NormArgs& a, hipStream_t s) { return pick_element(a, s, false); }
size_t norm_workspace_bytes(int width, int cus) { return (size_t)kParts * 2 * (size_t)width * sizeof(float); }

}  // namespace vkfx
