// linear_step.hip -- linear attention token by token: the recurrence itself.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "sequence.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

constexpr int kColumns = 16;             // state columns of a block
constexpr int kRowGroups = 16;           // threads along the rows of a column
constexpr int kRowsMost = 256 / kRowGroups;

// A block holds kColumns columns of one sequence's and head's state, a thread
// one column of every kRowGroups-th row, and walks the tokens.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_recurrent(const ScanArgs s, const float* __restrict__ powers) {
    __shared__ float part[kRowGroups][kColumns];
    const int h = blockIdx.y, b = blockIdx.z;
    const int col = threadIdx.x % kColumns, row0 = threadIdx.x / kColumns;
    const int c = blockIdx.x * kColumns + col;
    const bool live = c < s.dv;
    long long n = s.tokens;
    if (s.lengths) {
        const long long l = s.lengths[b];
        n = l < 0 ? 0 : l < n ? l : n;
    }
    // the decay in two parts: its rounding to 32 bits would grow with the
    // tokens that a long memory spans
    const float decay = powers[(long long)h * kDecayPowers + 1];
    const float decay_low = powers[(long long)h * kDecayPowers + kDecayPowers - 1];
    const long long st = ((long long)b * s.heads + h) * s.dk * s.dv;
    float x[kRowsMost];
#pragma unroll
    for (int k = 0; k < kRowsMost; ++k) {
        const int r = row0 + k * kRowGroups;
        x[k] = live && r < s.dk && s.state_in ? s.state_in[st + (long long)r * s.state_row + (long long)c * s.state_col] : 0.f;
    }
    const T* A = (const T*)s.a.p + b * s.a.batch + (h / s.a.group) * s.a.head;
    const T* B = (const T*)s.b.p + b * s.b.batch + (h / s.b.group) * s.b.head;
    const T* C = (const T*)s.c.p + b * s.c.batch + (h / s.c.group) * s.c.head;
    const long long ob = b * s.out_batch + h * s.out_head;
    for (long long i = 0; i < s.tokens; ++i) {
        const bool inside = i < n;
        const long long t = s.reverse && inside ? n - 1 - i : i;
        float o = 0.f;
        if (inside) {
            const float cv = live ? (float)C[t * s.c.token + c] * s.scale_update : 0.f;
#pragma unroll
            for (int k = 0; k < kRowsMost; ++k) {
                const int r = row0 + k * kRowGroups;
                if (r < s.dk) {
                    if (!s.reverse) x[k] = fmaf(x[k], decay, x[k] * decay_low);
                    x[k] = fmaf((float)B[t * s.b.token + r], cv, x[k]);
                    o = fmaf((float)A[t * s.a.token + r], x[k], o);
                    if (s.reverse) x[k] = fmaf(x[k], decay, x[k] * decay_low);
                }
            }
        }
        __syncthreads();
        part[row0][col] = o;
        __syncthreads();
        if (row0 == 0 && live) {
            float sum = 0.f;
            for (int g = 0; g < kRowGroups; ++g) sum += part[g][col];
            sum *= s.scale_in;
            const long long at = ob + t * s.out_token + c;
            if (s.out_f32) ((float*)s.out)[at] = sum;
            else ((T*)s.out)[at] = (T)sum;
        }
    }
    if (s.state_out)
#pragma unroll
        for (int k = 0; k < kRowsMost; ++k) {
            const int r = row0 + k * kRowGroups;
            if (live && r < s.dk) s.state_out[st + (long long)r * s.state_row + (long long)c * s.state_col] = x[k];
        }
}

}  // namespace

int launch_scan_recurrent(int element, const ScanArgs* scans, int count, const float* powers, hipStream_t s) {
    for (int i = 0; i < count; ++i) {
        const ScanArgs& a = scans[i];
        const dim3 grid((unsigned)((a.dv + kColumns - 1) / kColumns), (unsigned)a.heads, (unsigned)a.batch);
        if (element == VKFX_ELEMENT_F32) hipLaunchKernelGGL(k_scan_recurrent<float>, grid, dim3(256), 0, s, a, powers);
        else if (element == VKFX_ELEMENT_F16) hipLaunchKernelGGL(k_scan_recurrent<_Float16>, grid, dim3(256), 0, s, a, powers);
        else hipLaunchKernelGGL(k_scan_recurrent<__bf16>, grid, dim3(256), 0, s, a, powers);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return (int)hipSuccess;
}

}  // namespace vkfx
