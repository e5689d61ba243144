// linear_step.hip -- linear attention of one token of each sequence, or a few:
// the recurrence itself.
//
// Bound by memory: the state is read and written once, 8 dk dv bytes a head
// against 4 dk dv operations a token. A block holds CS columns of one head's
// state in its registers, four neighbours a lane and rows a fixed distance
// apart, and asks for all of them before it waits for any. Sums over the rows
// go through the lanes of a wave, then through LDS.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "sequence.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// CS columns a block, up to NR rows a thread. PACKED: a state's columns are
// neighbours in memory (they are not where a gradient reads its transpose).
// WHOLE: each thread has its NR rows.
template <typename T, int CS, int NR, bool PACKED, bool WHOLE>
__global__ __launch_bounds__(256) void k_step(const ScanArgs s, const float* __restrict__ powers) {
    constexpr int LX = CS / 4, RY = 256 / LX;  // lanes along a row, rows of the block
    __shared__ float la[kStepTokens][256], lb[kStepTokens][256], lc[kStepTokens][CS];
    __shared__ float part[kStepTokens][4][CS];
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int row0 = tid / LX, x0 = tid % LX * 4;
    const int col0 = blockIdx.x * CS, col = col0 + x0;
    int n = (int)s.tokens;
    if (s.lengths) n = s.lengths[b] < 0 ? 0 : s.lengths[b] < n ? s.lengths[b] : n;
    const long long st = ((long long)b * s.heads + h) * s.dk * s.dv;

    // Rows past the last read the last one again, for nothing: every load is on
    // its way before the first is waited for. Then they are zeros.
    f32x4 X[NR];
    const bool four = PACKED && col + 4 <= s.dv;
    if (!s.state_in) {
#pragma unroll
        for (int k = 0; k < NR; ++k) X[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    } else if (four) {
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int r = row0 + k * RY < s.dk ? row0 + k * RY : s.dk - 1;
            X[k] = *(const f32x4_any*)(s.state_in + st + (long long)r * s.state_row + col);
        }
    } else {
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int r = row0 + k * RY < s.dk ? row0 + k * RY : s.dk - 1;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                X[k][e] = col + e < s.dv ? s.state_in[st + (long long)r * s.state_row + (long long)(col + e) * s.state_col] : 0.f;
        }
    }
    // the tokens' rows, in the order of the scan
    const T* A = (const T*)s.a.p + b * s.a.batch + (h / s.a.group) * s.a.head;
    const T* B = (const T*)s.b.p + b * s.b.batch + (h / s.b.group) * s.b.head;
    const T* C = (const T*)s.c.p + b * s.c.batch + (h / s.c.group) * s.c.head;
    for (int i = 0; i < n; ++i) {
        const long long t = s.reverse ? n - 1 - i : i;
        la[i][tid] = tid < s.dk ? (float)A[t * s.a.token + tid] : 0.f;
        lb[i][tid] = tid < s.dk ? (float)B[t * s.b.token + tid] : 0.f;
        if (tid < CS) lc[i][tid] = col0 + tid < s.dv ? (float)C[t * s.c.token + col0 + tid] * s.scale_update : 0.f;
    }
    if constexpr (!WHOLE)
#pragma unroll
        for (int k = 0; k < NR; ++k)
            if (row0 + k * RY >= s.dk) X[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the decay in two parts, so that its rounding does not grow token by token
    const float decay = powers[(long long)h * kDecayPowers + kDecayHigh];
    const float decay_low = powers[(long long)h * kDecayPowers + kDecayLow];
    __syncthreads();
    // MASKED: rows past the last are left out; otherwise they meet zeros, which a value that is infinite would not survive.
    const auto advance = [&](int i, f32x4 c, f32x4& o, auto masked) {
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int r = row0 + k * RY;
            const float av = la[i][r], bv = lb[i][r];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = X[k][e];
                if (!s.reverse) x = fmaf(x, decay, x * decay_low);
                x = fmaf(bv, c[e], x);
                o[e] = !decltype(masked)::value || r < s.dk ? fmaf(av, x, o[e]) : o[e];
                if (s.reverse) x = fmaf(x, decay, x * decay_low);
                X[k][e] = decltype(masked)::value && r >= s.dk ? 0.f : x;
            }
        }
    };
    for (int i = 0; i < n; ++i) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        const f32x4 c = *(const f32x4*)&lc[i][x0];
        if (WHOLE || (c[0] * 0.f + c[1] * 0.f) + (c[2] * 0.f + c[3] * 0.f) == 0.f) advance(i, c, o, std::false_type{});
        else advance(i, c, o, std::true_type{});
#pragma unroll
        for (int d = LX; d < 64; d <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d);
        if ((tid & 63) < LX) *(f32x4*)&part[i][tid >> 6][x0] = o;
    }
    if (s.state_out && four) {
#pragma unroll
        for (int k = 0; k < NR; ++k)
            if (row0 + k * RY < s.dk) *(f32x4_any*)(s.state_out + st + (long long)(row0 + k * RY) * s.state_row + col) = X[k];
    } else if (s.state_out) {
#pragma unroll
        for (int k = 0; k < NR; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row0 + k * RY < s.dk && col + e < s.dv)
                    s.state_out[st + (long long)(row0 + k * RY) * s.state_row + (long long)(col + e) * s.state_col] = X[k][e];
    }
    __syncthreads();
    for (int j = tid; j < (int)s.tokens * CS; j += 256) {
        const int i = j / CS, c = j % CS;
        if (col0 + c >= s.dv) continue;
        const float y = i < n ? ((part[i][0][c] + part[i][1][c]) + (part[i][2][c] + part[i][3][c])) * s.scale_in : 0.f;
        const long long t = s.reverse && i < n ? n - 1 - i : i;
        const long long at = b * s.out_batch + t * s.out_token + h * s.out_head + col0 + c;
        if (s.out_f32) ((float*)s.out)[at] = y;
        else ((T*)s.out)[at] = (T)y;
    }
}

template <typename T, int CS, int NR>
void launch_as(const ScanArgs& a, const float* powers, hipStream_t s) {
    const dim3 grid((unsigned)((a.dv + CS - 1) / CS), (unsigned)a.heads, (unsigned)a.batch);
    const bool packed = a.state_col == 1, whole = a.dk == 256 * 4 / CS * NR;
    const auto kernel = packed ? (whole ? k_step<T, CS, NR, true, true> : k_step<T, CS, NR, true, false>)
                               : (whole ? k_step<T, CS, NR, false, true> : k_step<T, CS, NR, false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, powers);
}

// 64 columns a block; a fourth of that while those blocks would use less than an
// eighth of the CUs, where latency is a block's share of the state (4 heads of
// 256 x 256, 16 blocks of 64: 5.0 us, 4.2 with 16 columns; 32 blocks: 5.1 and 5.2;
// 16 heads of 128 x 128, 2 sequences, 64 blocks: 4.2 and 5.0, 32 sequences: 13.4
// and 23.6).
template <typename T>
void launch_element(const ScanArgs& a, const float* powers, int cus, hipStream_t s) {
    const long long blocks = (long long)a.batch * a.heads * ((a.dv + 63) / 64);
    if (blocks >= cus / 8) {
        if (a.dk <= 64) launch_as<T, 64, 4>(a, powers, s);
        else if (a.dk <= 128) launch_as<T, 64, 8>(a, powers, s);
        else launch_as<T, 64, 16>(a, powers, s);
    } else {
        if (a.dk <= 128) launch_as<T, 16, 2>(a, powers, s);
        else launch_as<T, 16, 4>(a, powers, s);
    }
}

}  // namespace

int launch_steps(int element, const ScanArgs* scans, int count, const float* powers, int cus, hipStream_t s) {
    for (int i = 0; i < count; ++i) {
        if (element == VKFX_ELEMENT_F32) launch_element<float>(scans[i], powers, cus, s);
        else if (element == VKFX_ELEMENT_F16) launch_element<_Float16>(scans[i], powers, cus, s);
        else launch_element<__bf16>(scans[i], powers, cus, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return (int)hipSuccess;
}

}  // namespace vkfx
