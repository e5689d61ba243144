// rotary.hip -- heads turned by their positions, with a norm of each in front
// where it is wanted, and the gradients of both.
//
// A pair (u1, u2) at position p turns by p f: (u1 c - u2 s, u1 s + u2 c); its
// gradient turns back, by -p f. f is kept as 64 bits of a turn, so p f is one
// product that wraps where an angle does, and its first bits are its quadrant:
// no position is too far. With the norm, n = x rstd, u = n weight:
//   du = the gradient turned back, g = du weight
//   dx = rstd (g - n mean(g n)),  dweight = sum du n
// over tokens and heads.
#include <algorithm>

#include "sequence.hpp"
#include "sequence_device.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

// Cosine and sine of 2^-64 `phase` turns, 1e-7 of each: the nearest quarter
// turn, then the series of what is left (to pi/4, the next term below 2^-32).
__device__ __forceinline__ void turn(uint64_t phase, float& c, float& s) {
    const unsigned quarter = ((unsigned)(phase >> 61) + 1) >> 1;
    const long long left = (long long)(phase - ((uint64_t)quarter << 62));
    const float t = fmaf((float)(unsigned)left, 0x1p-64f, (float)(int)(left >> 32) * 0x1p-32f);
    const float r = t * 6.283185307179586f, q = r * r;
    const float sn = r * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
    const float cs = fmaf(q, fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    c = quarter & 1 ? sn : cs;
    s = quarter & 1 ? cs : sn;
    if ((quarter + 1) & 2) c = -c;
    if (quarter & 2) s = -s;
}

__device__ __forceinline__ long long position(const RotaryArgs& a, long long b, long long t) {
    return a.positions ? a.positions[b * a.tokens + t] : a.starts ? a.starts[b] + t : t;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// A wave a row, up to 4 elements a lane, 64 apart. The block's sums of du n go
// to the workspace: row blockIdx.x of half blockIdx.y.
template <typename T, typename W, bool NORM, bool BACK>
__global__ __launch_bounds__(256) void k_rotary(const RotaryArgs a) {
    const RotaryRows& h = a.rows[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long rows = a.all * h.heads, stride = (long long)gridDim.x * 4;
    double sums[4] = {};
    for (long long r = (long long)blockIdx.x * 4 + wave; r < rows; r += stride) {
        const long long token = r / h.heads, b = token / a.tokens, t = token % a.tokens;
        const int head = (int)(r % h.heads);
        const T* x = (const T*)h.x.p + b * h.x.batch + t * h.x.token + head * h.x.head;
        T* out = (T*)h.out.p + b * h.out.batch + t * h.out.token + head * h.out.head;
        if (a.lengths && t >= a.lengths[b]) {
            for (int e = lane; e < a.dim; e += 64) out[e] = (T)0.f;
            continue;
        }
        const long long p = position(a, b, t);
        float v[4], w[4], c[4], s[4], n[4], other[4];
        float square = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = lane + 64 * j, half = a.turned / 2;
            v[j] = w[j] = c[j] = s[j] = n[j] = other[j] = 0.f;
            if (e >= a.dim) continue;
            v[j] = (float)x[e];
            w[j] = 1.f;
            if (NORM && h.weight) w[j] = (float)((const W*)h.weight)[e];
            c[j] = 1.f;
            if (e < a.turned) {
                const bool second = a.layout == VKFX_ROTARY_HALF ? e >= half : e & 1;
                const int pair = a.layout == VKFX_ROTARY_HALF ? e - second * half : e / 2;
                const int with = a.layout == VKFX_ROTARY_HALF ? (second ? pair : e + half) : e ^ 1;
                turn((uint64_t)p * a.turns[pair], c[j], s[j]);
                c[j] *= a.amplitude;
                s[j] *= second != BACK ? a.amplitude : -a.amplitude;
                other[j] = (float)x[with];
                if (NORM && !BACK && h.weight) other[j] *= (float)((const W*)h.weight)[with];
            }
            if constexpr (NORM && BACK) n[j] = (float)((const T*)h.in.p)[b * h.in.batch + t * h.in.token + head * h.in.head + e];
            square = NORM ? BACK ? fmaf(n[j], n[j], square) : fmaf(v[j], v[j], square) : 0.f;
        }
        float rstd = 1.f;
        if (NORM) {
            square = wave_sum(square);
            rstd = 1.f / sqrtf(square / (float)a.dim + a.epsilon);
            if (square == INFINITY) {  // squares past 32 bits: of 2^-68 of the row, beside which epsilon is nothing
                square = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float part = (BACK ? n[j] : v[j]) * 0x1p-68f;
                    square = fmaf(part, part, square);
                }
                rstd = 0x1p-68f / sqrtf(wave_sum(square) / (float)a.dim);
            }
        }
        if (!NORM || !BACK) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (lane + 64 * j < a.dim) out[lane + 64 * j] = (T)(fmaf(v[j] * w[j], c[j], other[j] * s[j]) * rstd);
            continue;
        }
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = fmaf(v[j], c[j], other[j] * s[j]);
            n[j] *= rstd;
            sums[j] += (double)(v[j] * n[j]);
            v[j] *= w[j];
            dot = fmaf(v[j], n[j], dot);
        }
        dot = wave_sum(dot) / (float)a.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) out[lane + 64 * j] = (T)((v[j] - n[j] * dot) * rstd);
    }
    if (!NORM || !BACK || !h.dweight) return;
    __shared__ double lds[4][256];
#pragma unroll
    for (int j = 0; j < 4; ++j) lds[wave][lane + 64 * j] = sums[j];
    __syncthreads();
    const int e = threadIdx.x;
    if (e < a.dim)
        a.partial[((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.dim + e] = (float)((lds[0][e] + lds[1][e]) + (lds[2][e] + lds[3][e]));
}

template <typename W>
__global__ __launch_bounds__(256) void k_rotary_weights(const RotaryArgs a, int parts) {
    const int e = threadIdx.x;
    W* to = (W*)a.rows[blockIdx.x].dweight;
    if (!to || e >= a.dim) return;
    double sum = 0.0;
    for (int i = 0; i < parts; ++i) sum += (double)a.partial[((long long)blockIdx.x * parts + i) * a.dim + e];
    to[e] = (W)(float)sum;
}

template <typename T, typename W, bool BACK>
int launch_as(const RotaryArgs& a, hipStream_t s) {
    const long long rows = a.all * std::max(a.rows[0].heads, a.rows[1].heads);
    const int blocks = (int)std::min((rows + 3) / 4, (long long)a.cus * 4);
    if (blocks) {
        if (a.norm) hipLaunchKernelGGL((k_rotary<T, W, true, BACK>), dim3(blocks, 2), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_rotary<T, W, false, BACK>), dim3(blocks, 2), dim3(256), 0, s, a);
    }
    if (BACK && (a.rows[0].dweight || a.rows[1].dweight))
        hipLaunchKernelGGL((k_rotary_weights<W>), dim3(2), dim3(256), 0, s, a, blocks);
    return (int)hipGetLastError();
}

template <typename T>
int pick(const RotaryArgs& a, hipStream_t s, bool back) {
    if (a.weight_element == VKFX_ELEMENT_F32) return back ? launch_as<T, float, true>(a, s) : launch_as<T, float, false>(a, s);
    return back ? launch_as<T, T, true>(a, s) : launch_as<T, T, false>(a, s);
}

int pick_element(const RotaryArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return pick<float>(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return pick<_Float16>(a, s, back);
    return pick<__bf16>(a, s, back);
}

}  // namespace

int launch_rotary_forward(const RotaryArgs& a, hipStream_t s) { return pick_element(a, s, false); }
int launch_rotary_backward(const RotaryArgs& a, hipStream_t s) { return pick_element(a, s, true); }
size_t rotary_workspace_bytes(int dim, int cus) { return (size_t)cus * 4 * 2 * (size_t)dim * sizeof(float); }

}  // namespace vkfx
